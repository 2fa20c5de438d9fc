"""The stand-alone operators on the GPU against their 64-bit statements (oracle/ops_ref.py).

Tolerances are elementwise and come from the statements: every rounding to bf16 moves a value by at most half a step
(2^-8 of it), a product of n terms summed in fp32 by at most n 2^-24 of the sum of absolute terms."""
import numpy as np
import pytest
import torch

from bidiff import ops
from oracle import ops_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def within(got, want, tol, what):
    got = got.detach().double()
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - want).abs() - tol
    assert float(over.max()) <= 1e-30, f"{what}: off by {float((got - want).abs().max()):.3g}, {float(over.max()):.3g} more than allowed"


# ------------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize("B,L,Hq,Hk,D,rd,inter,dt,how", [
    (1, 1, 1, 1, 32, 32, False, BF, "plain"), (2, 7, 3, 3, 64, 64, True, BF, "qkv"), (3, 5, 4, 2, 48, 24, False, BF, "qkv"),
    (2, 33, 5, 1, 128, 64, False, BF, "qkv"), (2, 33, 5, 1, 128, 64, True, torch.float32, "qkv"), (1, 9, 2, 2, 10, 6, True, BF, "plain"),
    (1, 9, 2, 2, 10, 6, False, torch.float32, "plain"), (2, 3, 2, 2, 80, 80, False, torch.float32, "qkv"), (4, 2, 12, 12, 64, 64, False, BF, "odd"),
    (2, 700, 40, 40, 64, 64, False, BF, "qkv"), (1, 6000, 16, 16, 128, 128, True, BF, "plain"), (2, 17, 3, 3, 64, 48, False, BF, "transposed"),
])
@pytest.mark.parametrize("given", [False, True])
def test_rotary_matches_the_formula(gpu_device, B, L, Hq, Hk, D, rd, inter, dt, how, given):
    dev, g = gpu_device, gen(gpu_device, B * L + D)
    n = max(L, 50)
    table = ops.rotary_table(rd, n, device=dev)

    def make(H):
        if how == "plain":
            return torch.randn(B, L, H, D, generator=g, device=dev).to(dt)
        if how == "transposed":      # [B, H, L, D] storage
            return torch.randn(B, H, L, D, generator=g, device=dev).to(dt).transpose(1, 2)
        x = torch.randn(B, L, H * D + (3 if how == "odd" else 16), generator=g, device=dev).to(dt)
        return x[..., 1 if how == "odd" else 8:][..., :H * D].unflatten(-1, (H, D))
    q, k = make(Hq).requires_grad_(True), make(Hk).requires_grad_(True)
    pos = torch.randint(0, n, (B, L), generator=g, device=dev) if given else None
    at = torch.arange(L, device=dev).expand(B, L) if pos is None else pos
    step = R.U if dt == BF else R.F

    def check(got, x, inverse, what):
        want = R.rotary(x.detach(), table, at, inter, inverse)
        terms = x.detach().double().abs()
        pair = R.rotary(terms, table.abs() * torch.tensor([1.0, -1.0], device=dev), at, inter)[..., :rd].abs()
        other = torch.cat([torch.maximum(pair, R.rotary(terms, table.abs(), at, inter)[..., :rd].abs()), terms[..., rd:]], -1)
        within(got, want, step * 1.01 * want.abs() + 4 * R.F * other, what)
        assert torch.equal(got[..., rd:], x.detach()[..., rd:])
    yq, yk = ops.rotary(q, k, table, pos, interleaved=inter)
    check(yq.detach(), q, False, "q")
    check(yk.detach(), k, False, "k")
    dq, dk = torch.randn_like(yq), torch.randn_like(yk)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    check(gq, dq, True, "dq")
    check(gk, dk, True, "dk")
    one, none = ops.rotary(q, None, table, pos, interleaved=inter)
    assert none is None and torch.equal(one, yq)
    (only,) = torch.autograd.grad(ops.rotary(q, k, table, pos, interleaved=inter)[1], (k,), (dk,))
    assert torch.equal(only, gk)
    with torch.no_grad():
        base = q.detach().clone(memory_format=torch.preserve_format)
        assert ops.rotary_(base, None, table, pos, interleaved=inter)[0] is base
        assert torch.equal(base, yq)


def test_rotary_rows_positions_outside_and_shared_positions(gpu_device):
    dev = gpu_device
    table = ops.rotary_table(16, 10, device=dev)
    x = torch.randn(6, 2, 32, device=dev)
    pos = torch.tensor([0, 9, 10, -1, 3, 2 ** 40], device=dev)
    y, _ = ops.rotary(x, None, table, pos)
    bad = torch.tensor([False, False, True, True, False, True], device=dev)
    assert bool(torch.isnan(y[bad][..., :16]).all()) and bool(torch.isfinite(y[~bad]).all()) and torch.equal(y[..., 16:], x[..., 16:])
    b = torch.randn(3, 4, 2, 32, device=dev).bfloat16()
    shared = torch.tensor([4, 1, 1, 8], device=dev)
    assert torch.equal(ops.rotary(b, None, table, shared)[0], ops.rotary(b, None, table, shared.expand(3, 4).contiguous())[0])
    assert torch.equal(ops.rotary(b, None, table, shared.expand(3, 4))[0], ops.rotary(b, None, table, shared)[0])
    far = ops.rotary_table(64, 131072, device=dev)          # a far position keeps fp32 accuracy
    z = torch.randn(1, 1, 1, 64, device=dev)
    at = torch.tensor([131071], device=dev)
    want = R.rotary(z, far, at[None], False)
    assert (ops.rotary(z, None, far, at)[0] - want).abs().max() < 4 * R.F * z.abs().max() * 2
    e, none = ops.rotary(b[:, :0], None, table)
    assert e.shape == (3, 0, 2, 32)


# ------------------------------------------------------------------------------------------------ differential attention
def attention_case(dev, B, Lq, Lk, H, Hkv, D, mask, lam, seed=0, scale_in=1.0, layout="plain"):
    g = gen(dev, seed + 1000 * B + Lq + 7 * Lk + H)
    rnd = lambda *s: (torch.randn(*s, generator=g, device=dev) * scale_in).to(BF)  # noqa: E731
    if layout == "qkv":            # one projection's output: q | k | v of a token side by side
        assert Lq == Lk
        x = rnd(B, Lq, 2 * H * D + 4 * Hkv * D)
        q, k, v = x.split([2 * H * D, 2 * Hkv * D, 2 * Hkv * D], -1)
        q, k, v = q.unflatten(-1, (2 * H, D)), k.unflatten(-1, (2 * Hkv, D)), v.unflatten(-1, (Hkv, 2 * D))
    elif layout == "heads":        # [B, heads, rows, D] storage
        q, k, v = (rnd(B, h, n, w).transpose(1, 2) for h, n, w in ((2 * H, Lq, D), (2 * Hkv, Lk, D), (Hkv, Lk, 2 * D)))
    elif layout == "odd":          # rows the kernels cannot read in 16-byte pieces: copied
        q, k, v = (rnd(B, n, h, w + 1)[..., 1:] for n, h, w in ((Lq, 2 * H, D), (Lk, 2 * Hkv, D), (Lk, Hkv, 2 * D)))
    else:
        q, k, v = rnd(B, Lq, 2 * H, D), rnd(B, Lk, 2 * Hkv, D), rnd(B, Lk, Hkv, 2 * D)
    lam = {"token": lambda: torch.rand(B, Lq, H, generator=g, device=dev).to(BF), "head": lambda: torch.rand(H, generator=g, device=dev),
           "row": lambda: torch.rand(B, Lq, 1, generator=g, device=dev), "one": lambda: torch.tensor(0.4, device=dev),
           "negative": lambda: -torch.rand(1, 1, H, generator=g, device=dev).to(BF), "batch": lambda: torch.rand(B, 1, H, generator=g, device=dev)}[lam]()
    m = None
    if mask == "tail":
        n = torch.randint(1, Lk + 1, (B,), generator=g, device=dev)
        m = torch.arange(Lk, device=dev)[None] < n[:, None]
    elif mask == "holes":
        m = torch.rand(B, Lk, generator=g, device=dev) < 0.5
    elif mask == "empty":
        m = torch.rand(B, Lk, generator=g, device=dev) < 0.5
        m[0] = False
    dout = rnd(B, Lq, H, 2 * D)
    return q, k, v, lam, m, dout


def reference(q, k, v, lam, m, dout, H):
    B, Lq, Lk = q.shape[0], q.shape[1], k.shape[1]
    full = lam.expand(B, Lq, H)
    spans = [(slice(b * Lq, (b + 1) * Lq), slice(b * Lk, (b + 1) * Lk)) for b in range(B)]
    seen = torch.ones(B * Lk, dtype=torch.bool, device=q.device) if m is None else m.reshape(-1) != 0
    flat = lambda x: None if x is None else x.detach().reshape(-1, *x.shape[2:])  # noqa: E731
    r = R.differential_attention(flat(q), flat(k), flat(v), flat(full), spans, seen, B * Lq, B * Lk, flat(dout), tol=True)
    return r


def lam_gradient(r, lam, lead, H):
    """(value, tolerance) of the gradient in lam's shape: sums over the axes it was broadcast along."""
    full, tol = r["dlam"].view(*lead, H), r["dlam_tol"].view(*lead, H)
    shape = (1,) * (3 - lam.dim()) + tuple(lam.shape)
    n = full.numel() / max(1, lam.numel())
    dims = [i for i in range(3) if shape[i] == 1 and full.shape[i] > 1]
    absolute = full.abs()
    for d in dims:
        full, tol, absolute = full.sum(d, keepdim=True), tol.sum(d, keepdim=True), absolute.sum(d, keepdim=True)
    step = R.U if lam.dtype == BF else R.F
    return full.reshape(lam.shape), (tol + absolute * (n + 8) * R.F + 1.01 * step * full.abs()).reshape(lam.shape)


SHAPES = [
    # B, Lq, Lk, H, Hkv, D, mask, lam, layout
    (1, 1, 1, 1, 1, 32, None, "token", "plain"), (2, 1, 2, 1, 1, 64, None, "head", "plain"), (1, 3, 65, 2, 1, 128, "holes", "row", "plain"),
    (2, 16, 16, 2, 2, 32, "empty", "token", "qkv"), (3, 17, 63, 2, 2, 64, "tail", "one", "plain"), (2, 64, 64, 3, 3, 64, "tail", "token", "qkv"),
    (2, 65, 64, 4, 2, 32, "holes", "negative", "heads"), (1, 127, 129, 2, 2, 64, None, "token", "odd"), (2, 128, 128, 3, 3, 64, "tail", "token", "qkv"),
    (1, 128, 128, 1, 1, 128, None, "token", "qkv"), (1, 129, 130, 4, 1, 128, "holes", "head", "plain"), (2, 200, 333, 2, 2, 64, "empty", "batch", "heads"),
    (1, 513, 511, 2, 1, 32, "tail", "token", "plain"), (1, 300, 700, 2, 2, 128, "holes", "token", "plain"), (5, 2, 700, 6, 3, 64, "tail", "token", "plain"),
    (1, 1, 3000, 8, 2, 64, "holes", "head", "plain"), (1, 4, 2500, 4, 1, 128, None, "token", "plain"), (1, 1, 5000, 1, 1, 32, "tail", "one", "plain"),
]


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,mask,lam,layout", SHAPES)
def test_differential_attention_forward_and_gradients(gpu_device, B, Lq, Lk, H, Hkv, D, mask, lam, layout):
    dev = gpu_device
    q, k, v, lam, m, dout = attention_case(dev, B, Lq, Lk, H, Hkv, D, mask, lam, layout=layout)
    r = reference(q, k, v, lam, m, dout, H)
    plain = ops.differential_attention(q, k, v, lam, key_mask=m)
    within(plain, r["out"].view(B, Lq, H, 2 * D), r["out_tol"].view(B, Lq, H, 2 * D), "out")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    out = ops.differential_attention(*leaves, key_mask=None if m is None else m.long())
    within(out.detach(), r["out"].view(out.shape), r["out_tol"].view(out.shape), "out (training)")
    grads = torch.autograd.grad(out, leaves, dout)
    for name, x, leaf in zip(("dq", "dk", "dv"), grads, leaves):
        assert x.dtype == BF and x.shape == leaf.shape
        within(x, r[name].view(x.shape), r[name + "_tol"].view(x.shape), name)
    want, tol = lam_gradient(r, lam, (B, Lq), H)
    assert grads[3].dtype == lam.dtype
    within(grads[3], want, tol, "dlam")
    again = torch.autograd.grad(ops.differential_attention(*leaves, key_mask=m), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))            # equal calls, equal bits
    if m is not None:      # masked places: nothing they hold reaches anything, their gradients are exact zeros
        for x in (grads[1], grads[2]):
            assert not bool(x[~m].any())
        empty = ~m.any(1)
        assert not bool(plain[empty].any()) and not bool(grads[0][empty].any())
        bad = [t.detach().clone() for t in (k, v)]
        for t, junk in zip(bad, (float("nan"), float("inf"))):
            t[~m] = junk
        bad = [t.requires_grad_(True) for t in bad]
        out2 = ops.differential_attention(leaves[0], *bad, leaves[3], key_mask=m)
        assert torch.equal(out2, out)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out2, (leaves[0], *bad, leaves[3]), dout), grads))


@pytest.mark.parametrize("lens,total,H,Hkv,D,masked", [
    ([1], 1, 1, 1, 64, False), ([0, 5, 0, 1, 64, 0], 70, 2, 2, 32, False), ([65, 128, 3], 256, 3, 3, 64, True), ([300, 0, 129, 7], 436, 2, 1, 128, False),
    ([0, 0], 6, 2, 2, 64, False), ([200, 190, 1, 77], 500, 4, 4, 32, True), ([31, 64, 2, 0, 17], 128, 6, 3, 64, False),
])
def test_differential_attention_packed_rows(gpu_device, lens, total, H, Hkv, D, masked):
    dev = gpu_device
    g = gen(dev, total + D)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)  # noqa: E731
    q, k, v, dout = rnd(total, 2 * H, D), rnd(total, 2 * Hkv, D), rnd(total, Hkv, 2 * D), rnd(total, H, 2 * D)
    lam = torch.rand(total, H, generator=g, device=dev).to(BF)
    cu = np.concatenate([[0], np.cumsum(lens)])
    cut = torch.tensor(cu, dtype=torch.int32, device=dev)
    longest = max(max(lens), 1)
    spans = [(slice(a, b), slice(a, b)) for a, b in zip(cu[:-1].tolist(), cu[1:].tolist())]
    seen, m = torch.ones(total, dtype=torch.bool, device=dev), None
    if masked:
        m = torch.rand(len(lens), longest, generator=g, device=dev) < 0.7
        for b, (a, e) in enumerate(zip(cu[:-1], cu[1:])):
            seen[a:e] = m[b, :e - a]
    r = R.differential_attention(q, k, v, lam, spans, seen, total, total, dout, tol=True)
    leaves = [t.requires_grad_(True) for t in (q, k, v, lam)]
    out = ops.differential_attention(*leaves, key_mask=m, cu_seqlens=cut, max_seqlen=longest)
    within(out.detach(), r["out"], r["out_tol"], "out")
    grads = torch.autograd.grad(out, leaves, dout)
    for name, x in zip(("dq", "dk", "dv"), grads):
        within(x, r[name], r[name + "_tol"], name)
    within(grads[3], r["dlam"], r["dlam_tol"] + 1.01 * R.U * r["dlam"].abs(), "dlam")
    for x in (out, *grads):                                                # rows behind the last sequence
        assert not bool(x[cu[-1]:].any())
    if sum(lens):
        assert torch.equal(ops.differential_attention(*[t.detach() for t in leaves], key_mask=m, cu_seqlens=cut.long()), out)
        head = torch.rand(H, generator=g, device=dev).requires_grad_(True)     # a weight per head: its gradient sums over rows
        full = head.detach().expand(total, H)
        r2 = R.differential_attention(q, k, v, full, spans, seen, total, total, dout, tol=True)
        (dh,) = torch.autograd.grad(ops.differential_attention(q, k, v, head, key_mask=m, cu_seqlens=cut, max_seqlen=longest), (head,), dout)
        within(dh, r2["dlam"].sum(0), r2["dlam_tol"].sum(0) + r2["dlam"].abs().sum(0) * (total + 8) * R.F + R.F * r2["dlam"].sum(0).abs(), "dlam by head")


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [
    (1, 1, 1, 1, 1, 64), (3, 5, 1, 4, 2, 32), (4, 70, 1, 2, 1, 128), (2, 9, 40, 2, 2, 64), (3, 129, 128, 3, 3, 64), (2, 20, 200, 4, 1, 64),
    (2, 33, 300, 2, 2, 32), (2, 300, 150, 2, 1, 128), (2, 17, 1100, 2, 2, 128),
])
def test_differential_attention_one_key_seen(gpu_device, B, Lq, Lk, H, Hkv, D):
    """One key has weight 1 whatever its score: out = (1 - lam) v, and q and k have a gradient of exactly zero."""
    dev = gpu_device
    q, k, v, lam, _, dout = attention_case(dev, B, Lq, Lk, H, Hkv, D, None, "token")
    m = torch.zeros(B, Lk, dtype=torch.bool, device=dev)
    m[torch.arange(B), torch.arange(B) * 37 % Lk] = True
    r = reference(q, k, v, lam, m, dout, H)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    for mask in (m, None) if Lk == 1 else (m,):
        out = ops.differential_attention(*leaves, key_mask=mask)
        within(out.detach(), r["out"].view(out.shape), r["out_tol"].view(out.shape), "out")
        dq, dk, dv, dlam = torch.autograd.grad(out, leaves, dout)
        assert not bool(dq.any()) and not bool(dk.any())
        within(dv, r["dv"].view(dv.shape), r["dv_tol"].view(dv.shape), "dv")
        want, tol = lam_gradient(r, lam, (B, Lq), H)
        within(dlam, want, tol, "dlam")
    if Lk > 1:                                             # a second key for the last entry: its gradients are back, the others' stay zero
        m[-1, (B * 37 - 36) % Lk] = True
        r = reference(q, k, v, lam, m, dout, H)
        dq, dk = torch.autograd.grad(ops.differential_attention(*leaves, key_mask=m), leaves[:2], dout)
        assert not bool(dq[:-1].any()) and not bool(dk[:-1].any()) and bool(dq[-1].any()) and bool(dk[-1].any())
        within(dq, r["dq"].view(dq.shape), r["dq_tol"].view(dq.shape), "dq")
        within(dk, r["dk"].view(dk.shape), r["dk_tol"].view(dk.shape), "dk")


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [(2, 60, 300, 2, 1, 32), (1, 130, 513, 2, 2, 64), (1, 40, 1100, 1, 1, 128), (2, 60, 120, 2, 1, 32), (1, 40, 400, 2, 2, 64)])
def test_differential_attention_weight_gradient_keeps_fp32(gpu_device, B, Lq, Lk, H, Hkv, D):
    """Every value row holds x in one column: a row's dlam is -x dout of that column, with no error of weights in bf16
    (about 1e-4 here). Relative: both sums over the keys Lk steps of 2^-24, the scores' dot products D steps of their
    absolute sum in each pass, the exponents a step of their size."""
    dev = gpu_device
    q, k, _, _, _, dout = attention_case(dev, B, Lq, Lk, H, Hkv, D, None, "token")
    v = torch.zeros(B, Lk, Hkv, 2 * D, dtype=BF, device=dev)
    v[..., 5] = 1.5
    lam = torch.full((B, Lq, H), 0.5, device=dev, requires_grad=True)
    out = ops.differential_attention(q.requires_grad_(True), k, v, lam)
    (dlam,) = torch.autograd.grad(out, (lam,), dout)
    want = -1.5 * dout[..., 5].double()
    absolute = float((q.detach().float().norm(dim=-1).max() * k.float().norm(dim=-1).max()).item()) / D ** 0.5
    rel = R.F * (2 * Lk + 2 * D * absolute + 8 * absolute + 16)
    within(dlam, want, rel * want.abs(), "dlam")


@pytest.mark.parametrize("lens,D", [([1], 32), ([1] * 9, 64), ([1, 0, 1, 1], 128), ([1, 2, 1, 70, 1], 64)])
def test_differential_attention_packed_rows_of_one_token(gpu_device, lens, D):
    dev, total, H, Hkv = gpu_device, sum(lens) + 2, 4, 2
    g = gen(dev, total + D)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF)  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (rnd(total, 2 * H, D), rnd(total, 2 * Hkv, D), rnd(total, Hkv, 2 * D), rnd(total, H))]
    cu = torch.tensor([0, *np.cumsum(lens)], dtype=torch.int32, device=dev)
    out = ops.differential_attention(*leaves, cu_seqlens=cu)
    dq, dk, dv, _ = torch.autograd.grad(out, leaves, rnd(total, H, 2 * D))
    alone = torch.zeros(total, dtype=torch.bool, device=dev)
    for n, at in zip(lens, cu.tolist()):
        alone[at:at + n] = n == 1
    assert not bool(dq[alone].any()) and not bool(dk[alone].any()) and bool(dv[alone].any())
    seen = ~alone & (torch.arange(total, device=dev) < cu[-1])
    assert bool((dq[seen].flatten(1) != 0).any(1).all()) and bool((dk[seen].flatten(1) != 0).any(1).all())


def test_differential_attention_packed_rows_longer_than_announced_are_nan(gpu_device):
    dev = gpu_device
    x = [torch.randn(20, h, w, device=dev).to(BF) for h, w in ((4, 32), (4, 32), (2, 64))]
    cu = torch.tensor([0, 4, 16, 20], dtype=torch.int32, device=dev)
    out = ops.differential_attention(*x, torch.tensor(0.3, device=dev), cu_seqlens=cu, max_seqlen=8)
    assert bool(torch.isnan(out[12:16]).all()) and bool(torch.isfinite(out[:12]).all()) and bool(torch.isfinite(out[16:]).all())


def test_differential_attention_packed_rows_of_no_sequence(gpu_device):
    """Zeros before the first and behind the last sequence; in a sequence longer than announced NaN from there on, in every
    gradient as well; the rows of the other sequences as if they were alone."""
    dev, g = gpu_device, gen(gpu_device, 21)
    x = [torch.randn(70, h, w, generator=g, device=dev).to(BF).requires_grad_(True) for h, w in ((4, 32), (4, 32), (2, 64))]
    lam = torch.rand(70, 2, generator=g, device=dev).requires_grad_(True)
    dout = torch.randn(70, 2, 64, generator=g, device=dev).to(BF)
    cu = torch.tensor([3, 9, 9, 40, 60], dtype=torch.int32, device=dev)
    out = ops.differential_attention(*x, lam, cu_seqlens=cu, max_seqlen=25)
    grads = torch.autograd.grad(out, (*x, lam), dout)
    for y in (out.detach(), *grads):
        assert not bool(y[:3].any()) and not bool(y[60:].any())
        assert bool(torch.isnan(y[34:40].float()).all()) and bool(torch.isfinite(y[:34].float()).all()) and bool(torch.isfinite(y[40:].float()).all())
    for a, b in ((3, 9), (40, 60)):
        one = [t.detach()[a:b].requires_grad_(True) for t in (*x, lam)]
        alone = ops.differential_attention(*one, cu_seqlens=torch.tensor([0, b - a], dtype=torch.int32, device=dev), max_seqlen=25)
        assert torch.equal(alone, out[a:b])
        assert all(torch.equal(s, t[a:b]) for s, t in zip(torch.autograd.grad(alone, one, dout[a:b]), grads))


def test_differential_attention_without_rows_or_keys(gpu_device):
    dev = gpu_device
    for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        t = [torch.zeros(B, n, h, w, dtype=BF, device=dev, requires_grad=True) for n, h, w in ((Lq, 4, 32), (Lk, 4, 32), (Lk, 2, 64))]
        lam = torch.zeros(2, device=dev, requires_grad=True)
        out = ops.differential_attention(*t, lam)
        assert out.shape == (B, Lq, 2, 64) and not bool(out.any())
        out.sum().backward()
        assert all(x.grad is not None and not bool(x.grad.any()) for x in (*t, lam))


def test_differential_attention_extreme_scores(gpu_device):
    """Scores far apart (one key takes all weight) and uniform attention with a common value (the gradients are small
    differences): both stay within the bounds."""
    dev = gpu_device
    for Lk in (100, 400):
        q, k, v, lam, m, dout = attention_case(dev, 1, 70, Lk, 2, 2, 64, None, "token", seed=9, scale_in=6.0)
        for scale_in, vv in ((1.0, v), (0.0, (v.float() * 0.1 + 5.0).to(BF))):
            qq = (q.float() * scale_in).to(BF)
            r = reference(qq, k, vv, lam, m, dout, 2)
            leaves = [t.detach().requires_grad_(True) for t in (qq, k, vv, lam)]
            out = ops.differential_attention(*leaves)
            within(out.detach(), r["out"].view(out.shape), r["out_tol"].view(out.shape), "out")
            for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)):
                within(x, r[name].view(x.shape), r[name + "_tol"].view(x.shape), name)


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,mask,lam", [
    (1, 40, 2100, 2, 2, 64, "holes", "token"), (2, 33, 2049, 4, 2, 64, "empty", "head"), (1, 70, 4200, 4, 1, 128, None, "token"), (1, 100, 3300, 2, 1, 32, "tail", "row"),
    (1, 16, 9000, 4, 1, 64, None, "token"), (1, 9, 1200, 6, 1, 128, "holes", "token"), (3, 5, 260, 3, 3, 32, "tail", "negative"), (1, 31, 2048, 1, 1, 64, "holes", "one"),
])
def test_differential_attention_split_over_keys(gpu_device, B, Lq, Lk, H, Hkv, D, mask, lam):
    """Workgroups of either size with their keys split, joined from few and from many splits; splits without a visible key."""
    q, k, v, lm, m, dout = attention_case(gpu_device, B, Lq, Lk, H, Hkv, D, mask, lam, seed=Lk)
    r = reference(q, k, v, lm, m, dout, H)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lm)]
    out = ops.differential_attention(*leaves, m)
    within(out.detach(), r["out"].view(out.shape), r["out_tol"].view(out.shape), "out")
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, dout)):
        within(x, r[name].view(x.shape), r[name + "_tol"].view(x.shape), name)
    with torch.no_grad():
        assert torch.equal(ops.differential_attention(*leaves, m), out)


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,mask", [
    (70, 65, 64, 2, 2, 64, "holes"), (44, 130, 520, 3, 3, 64, "tail"), (66, 129, 130, 2, 1, 128, "empty"), (33, 100, 1030, 4, 4, 128, None), (150, 40, 70, 4, 2, 32, "tail"),
    (70, 65, 140, 2, 2, 64, "holes"), (3, 70, 200, 2, 1, 64, "empty"), (80, 70, 129, 2, 2, 32, "empty"), (20, 128, 128, 6, 2, 64, "holes"),
])
def test_differential_attention_many_workgroups(gpu_device, B, Lq, Lk, H, Hkv, D, mask):
    """Enough queries for every CU: the larger workgroups of the query side's gradient, keys walked once and twice."""
    q, k, v, lm, m, dout = attention_case(gpu_device, B, Lq, Lk, H, Hkv, D, mask, "token", seed=B + D)
    r = reference(q, k, v, lm, m, dout, H)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lm)]
    out = ops.differential_attention(*leaves, m)
    within(out.detach(), r["out"].view(out.shape), r["out_tol"].view(out.shape), "out")
    grads = torch.autograd.grad(out, leaves, dout)
    for name, x in zip(("dq", "dk", "dv"), grads):
        within(x, r[name].view(x.shape), r[name + "_tol"].view(x.shape), name)
    want, tol = lam_gradient(r, lm, (B, Lq), H)
    within(grads[3], want, tol, "dlam")
    again = torch.autograd.grad(ops.differential_attention(*leaves, m), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("shape", [(), (1,), (3,), (1, 3), (70, 1), (70, 3), (1, 70, 1), (1, 1, 3), (150, 1, 1), (150, 1, 3), (150, 70, 1), (1, 70, 3), (1, 1, 1)])
def test_differential_attention_broadcast_weights(gpu_device, shape):
    """The gradient of a weight that is shared along any axes is the sum of the gradients it has where it is not."""
    dev, g = gpu_device, gen(gpu_device, 31)
    q, k, v = (torch.randn(150, 70, h, w, generator=g, device=dev).to(BF) for h, w in ((6, 32), (6, 32), (3, 64)))
    dout = torch.randn(150, 70, 3, 64, generator=g, device=dev).to(BF)
    lam = torch.rand(shape, generator=g, device=dev)
    full = lam.expand(150, 70, 3).contiguous().requires_grad_(True)
    (want,) = torch.autograd.grad(ops.differential_attention(q, k, v, full), (full,), dout)
    lam.requires_grad_(True)
    out = ops.differential_attention(q, k, v, lam)
    (got,) = torch.autograd.grad(out, (lam,), dout)
    assert got.shape == lam.shape and got.dtype == torch.float32
    dims = [d for d, n in enumerate((1,) * (3 - len(shape)) + tuple(shape)) if n == 1]
    total, size = (x.double().sum(dims, keepdim=True).reshape(shape) for x in (want, want.abs()))
    n = want.numel() // max(1, lam.numel())
    # n - 1 additions in fp32, every partial sum at most the sum of the sizes
    assert bool(((got.double() - total).abs() <= n * R.F * size).all())


def test_differential_attention_long_cache_offsets(gpu_device):
    """Keys whose byte offset passes 32 bits: rows of a buffer of more than 4 GiB, strided."""
    dev = gpu_device
    rows, stride = 4096, 600_000                       # 4096 rows of 1.2 MB: 4.9 GB
    buf = torch.empty(rows * stride, dtype=BF, device=dev)
    g = gen(dev, 77)
    k = buf.as_strided((1, rows, 2, 64), (rows * stride, stride, 64, 1))
    v = buf.as_strided((1, rows, 1, 128), (rows * stride, stride, 128, 1), 128)
    k.copy_(torch.randn(1, rows, 2, 64, generator=g, device=dev))
    v.copy_(torch.randn(1, rows, 1, 128, generator=g, device=dev))
    q = torch.randn(1, 3, 2, 64, generator=g, device=dev).to(BF)
    lam = torch.tensor(0.7, device=dev)
    a = ops.differential_attention(q, k, v, lam)
    b = ops.differential_attention(q, k.contiguous(), v.contiguous(), lam)
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ vocabulary head
@pytest.mark.parametrize("M,d,V,live,wdt", [
    (1, 64, 1, 1.0, BF), (1, 64, 2, 1.0, BF), (3, 128, 39, 0.7, BF), (64, 192, 63, 0.5, torch.float32), (65, 64, 64, 1.0, BF), (130, 384, 65, 0.5, BF),
    (257, 384, 803, 0.5, torch.float32), (1000, 320, 1025, 0.1, BF), (300, 2048, 130, 0.9, BF), (2049, 128, 5003, 0.5, BF), (40, 64, 70001, 0.5, BF),
    (9000, 64, 9001, 0.6, BF),
])
def test_linear_cross_entropy(gpu_device, M, d, V, live, wdt):
    dev, g = gpu_device, gen(gpu_device, M + d + V)
    h = torch.randn(M, d, generator=g, device=dev).to(BF)
    e = (torch.randn(V, d, generator=g, device=dev) * 2.0 / d ** 0.5).to(wdt)
    t = torch.randint(0, V, (M,), generator=g, device=dev)
    ind = torch.rand(M, generator=g, device=dev) < live
    ind[0] = True
    am = (torch.rand(M, generator=g, device=dev) < 0.8).long()
    am[0] = 1
    w = ind.float() * am.float()
    h[w == 0] = float("nan")                       # rows without weight are never read
    t[w == 0] = -100
    r = R.linear_cross_entropy(torch.where(w[:, None] > 0, h, torch.zeros_like(h)), e.to(BF), torch.where(w > 0, t, torch.zeros_like(t)), w, gout=0.25, tol=True)
    leaves = [h.requires_grad_(True), e.requires_grad_(True)]
    loss = ops.linear_cross_entropy(*leaves, t, ind, am)
    within(loss.detach(), r["loss"], r["loss_tol"], "loss")
    dh, de = torch.autograd.grad(loss / 4, leaves)
    assert dh.dtype == BF and de.dtype == wdt
    within(dh, r["dh"], r["dh_tol"], "dhidden")
    within(de, r["dw"], r["dw_tol"], "dweight")
    assert not bool(dh[w == 0].any())
    with torch.no_grad():
        assert torch.equal(ops.linear_cross_entropy(*leaves, t, ind, am), loss)
    again = torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, ind, am) / 4, leaves)
    assert torch.equal(again[0], dh) and torch.equal(again[1], de)


@pytest.mark.parametrize("M,d,V,live,wdt", [(5000, 1024, 65000, 0.3, BF), (9000, 256, 65000, 0.2, torch.float32)])
def test_linear_cross_entropy_in_pieces_of_the_vocabulary(gpu_device, M, d, V, live, wdt):
    """The largest tiles of every product, and a backward in several pieces of the vocabulary."""
    dev, g = gpu_device, gen(gpu_device, M + V)
    h = torch.randn(M, d, generator=g, device=dev).to(BF)
    e = (torch.randn(V, d, generator=g, device=dev) * 2.0 / d ** 0.5).to(wdt)
    t = torch.randint(0, V, (M,), generator=g, device=dev)
    ind = torch.rand(M, generator=g, device=dev) < live
    rows = ind.nonzero()[:, 0]
    r = R.linear_cross_entropy(h[rows], e.to(BF), t[rows], torch.ones(len(rows), device=dev), gout=1.0, tol=True)
    leaves = [h.requires_grad_(True), e.requires_grad_(True)]
    loss = ops.linear_cross_entropy(*leaves, t, ind)
    within(loss.detach(), r["loss"], r["loss_tol"], "loss")
    dh, de = torch.autograd.grad(loss, leaves)
    within(dh[rows], r["dh"], r["dh_tol"], "dhidden")
    within(de, r["dw"], r["dw_tol"], "dweight")
    assert not bool(dh[~ind].any())
    again = torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, ind), leaves)
    assert torch.equal(again[0], dh) and torch.equal(again[1], de)


def test_linear_cross_entropy_agrees_with_the_logits_form(gpu_device):
    """The same value as masked_cross_entropy on the product's logits, [B, L] shapes, fp32 hidden, without masks."""
    from bidiff.training.autograd import masked_cross_entropy
    dev, g = gpu_device, gen(gpu_device, 5)
    h = torch.randn(4, 33, 128, generator=g, device=dev).to(BF).float().requires_grad_(True)
    e = (torch.randn(71, 128, generator=g, device=dev) * 0.1).to(BF)
    t = torch.randint(0, 71, (4, 33), generator=g, device=dev)
    ind, am = torch.rand(4, 33, generator=g, device=dev) < 0.4, (torch.rand(4, 33, generator=g, device=dev) < 0.9).long()
    logits = (h.detach() @ e.float().t())
    for i, a in ((ind, am), (ind, None), (ind.to(torch.int32) * 256, am.int())):
        want = masked_cross_entropy(logits, t, i != 0, None if a is None else a.long())
        got = ops.linear_cross_entropy(h, e, t, i, a)
        assert abs(float(got - want)) < 1e-5 * max(1.0, float(want))
    both = ops.linear_cross_entropy(h, e, t)
    want = torch.nn.functional.cross_entropy(logits.view(-1, 71), t.view(-1))
    assert abs(float(both - want)) < 1e-5 * float(want)
    (dh,) = torch.autograd.grad(both, (h,))
    assert dh.dtype == torch.float32 and dh.shape == h.shape


def test_linear_cross_entropy_without_rows_and_with_bad_targets(gpu_device):
    dev = gpu_device
    h = torch.randn(70, 64, device=dev).to(BF).requires_grad_(True)
    e = torch.randn(9, 64, device=dev).to(BF).requires_grad_(True)
    t = torch.zeros(70, dtype=torch.long, device=dev)
    zero = ops.linear_cross_entropy(h, e, t, torch.zeros(70, dtype=torch.bool, device=dev))
    zero.backward()
    assert zero.item() == 0.0 and not bool(h.grad.any()) and not bool(e.grad.any())
    none = ops.linear_cross_entropy(h[:0], e, t[:0])
    none.backward()
    assert none.item() == 0.0
    for bad in (-1, 9, 2 ** 40):
        t2 = t.clone()
        t2[3] = bad
        assert bool(torch.isnan(ops.linear_cross_entropy(h, e, t2)))
        live = torch.ones(70, device=dev)
        live[3] = 0
        assert bool(torch.isfinite(ops.linear_cross_entropy(h, e, t2, live)))
