"""The 64-bit statements of the stand-alone operators against themselves: written gradients against central differences
and against autograd of an independent expression, on the CPU."""
import math

import numpy as np
import pytest
import torch

from oracle import ops_ref as R


def central(f, x, dy, eps=1e-6):
    """Directional derivatives of <f(x), dy> for every entry of x."""
    g = torch.zeros_like(x)
    flat, gf = x.view(-1), g.view(-1)
    for i in range(flat.numel()):
        keep = flat[i].item()
        flat[i] = keep + eps
        up = (f() * dy).sum()
        flat[i] = keep - eps
        down = (f() * dy).sum()
        flat[i] = keep
        gf[i] = (up - down) / (2 * eps)
    return g


@pytest.mark.parametrize("Hkv,share", [(1, 1), (1, 2), (2, 1)])
def test_differential_attention_gradients_against_differences(Hkv, share):
    g = torch.Generator().manual_seed(Hkv * 10 + share)
    Lq, Lk, H, D = 3, 5, Hkv * share, 4
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, lam, dout = rnd(Lq, 2 * H, D), rnd(Lk, 2 * Hkv, D), rnd(Lk, Hkv, 2 * D), rnd(Lq, H), rnd(Lq, H, 2 * D)
    seen = torch.tensor([True, True, False, True, True])
    call = lambda d=None: R.differential_attention(q, k, v, lam, [(slice(0, Lq), slice(0, Lk))], seen, Lq, Lk, d)  # noqa: E731
    r = call(dout)
    for name, x in (("dq", q), ("dk", k), ("dv", v), ("dlam", lam)):
        want = central(lambda: call()["out"], x, dout)
        assert (r[name] - want).abs().max() < 1e-7, name
    assert float(r["dk"][2].abs().max()) == 0.0 and float(r["dv"][2].abs().max()) == 0.0


def test_differential_attention_row_without_keys_and_garbage_behind_the_mask():
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 2, 4), (3, 2, 4), (3, 1, 8)))
    lam = torch.full((2, 1), 0.5, dtype=torch.float64)
    spans = [(slice(0, 2), slice(0, 3))]
    none = R.differential_attention(q, k, v, lam, spans, torch.zeros(3, dtype=torch.bool), 2, 3, torch.ones(2, 1, 8))
    assert all(float(x.abs().max()) == 0.0 for x in none.values())
    k[1], v[1] = math.nan, math.inf
    some = R.differential_attention(q, k, v, lam, spans, torch.tensor([True, False, True]), 2, 3, torch.ones(2, 1, 8))
    assert all(bool(torch.isfinite(x).all()) for x in some.values())


def test_linear_cross_entropy_gradients_against_differences():
    g = torch.Generator().manual_seed(4)
    M, d, V = 6, 5, 7
    h, e = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((M, d), (V, d)))
    t = torch.randint(0, V, (M,), generator=g)
    w = torch.tensor([1.0, 0.0, 1.0, 1.0, 0.0, 1.0], dtype=torch.float64)
    one = torch.tensor(1.7, dtype=torch.float64)
    r = R.linear_cross_entropy(h, e, t, w, gout=1.7)
    f = lambda: R.linear_cross_entropy(h, e, t, w)["loss"]  # noqa: E731
    assert (r["dh"] - central(f, h, one)).abs().max() < 1e-8
    assert (r["dw"] - central(f, e, one)).abs().max() < 1e-8
    want = torch.nn.functional.cross_entropy((h @ e.t())[w > 0], t[w > 0])
    assert abs(float(r["loss"] - want)) < 1e-12
    zero = R.linear_cross_entropy(h, e, t, torch.zeros(M))
    assert float(zero["loss"]) == 0.0 and float(zero["dh"].abs().max()) == 0.0


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_is_a_rotation_and_its_gradient_turns_back(interleaved):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 3, 2, 10, generator=g, dtype=torch.float64)
    ang = torch.rand(8, 3, generator=g, dtype=torch.float64) * 6
    table = torch.stack([ang.cos(), ang.sin()], -1)
    pos = torch.tensor([[0, 5, 7], [2, 2, 1]])
    y = R.rotary(x, table, pos, interleaved)
    assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[..., 6:], x[..., 6:])
    dy = torch.randn(*x.shape, generator=g, dtype=torch.float64)
    want = central(lambda: R.rotary(x, table, pos, interleaved), x, dy)
    assert (R.rotary(dy, table, pos, interleaved, inverse=True) - want).abs().max() < 1e-8
    assert torch.allclose(R.rotary(y, table, pos, interleaved, inverse=True), x)
    assert bool(torch.isnan(R.rotary(x, table, torch.full((2, 3), 8), interleaved)[..., :6]).all())


def test_rotary_table_rules_in_64_bits():
    """Entries against angles of their own: far positions keep the accuracy of their fp32 rounding (2^-24), linear
    stretching is the plain table at divided positions, ntk keeps the fastest pair and stretches the slowest by the
    factor, yarn keeps fast pairs, stretches slow ones and scales by 0.1 ln(factor) + 1."""
    from bidiff import ops
    n, dim = 200001, 16
    f = 10000.0 ** (-2.0 * np.arange(8) / dim)
    t = ops.rotary_table(dim, n).double().numpy()
    for pos in (0, 1, 4097, 200000):
        assert np.abs(t[pos, :, 0] - np.cos(pos * f)).max() < 1.01 * 2.0 ** -24 + 1e-10
        assert np.abs(t[pos, :, 1] - np.sin(pos * f)).max() < 1.01 * 2.0 ** -24 + 1e-10
    lin = ops.rotary_table(dim, 4001, scaling="linear", factor=4.0)
    assert torch.allclose(lin[::4], ops.rotary_table(dim, 1001), atol=1e-6)
    ntk = ops.rotary_table(dim, 3, scaling="ntk", factor=8.0).double().numpy()
    fn = np.arctan2(ntk[1, :, 1], ntk[1, :, 0])
    assert abs(fn[0] - f[0]) < 1e-6 and abs(fn[-1] * 8.0 / f[-1] - 1.0) < 1e-3
    ya = ops.rotary_table(64, 3, scaling="yarn", factor=4.0, original_positions=4096).double().numpy()
    fy, f64 = np.arctan2(ya[1, :, 1], ya[1, :, 0]), 10000.0 ** (-2.0 * np.arange(32) / 64)
    assert np.allclose(np.hypot(ya[1, :, 0], ya[1, :, 1]), 0.1 * math.log(4.0) + 1.0, atol=1e-6)
    assert abs(fy[0] - f64[0]) < 1e-6 and abs(fy[-1] / (f64[-1] / 4.0) - 1.0) < 1e-3
    assert np.all(fy <= f64 * (1 + 1e-6)) and np.all(fy >= f64 / 4.0 * (1 - 1e-3))
